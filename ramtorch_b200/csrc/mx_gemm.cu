// Products of microscaled operands on the fifth-generation tensor cores: the weight gradient from
// an 8-bit checkpoint, and the product of two MXFP4 matrices.
//
// Both compute the transposed output tile: the 128 lanes of the accumulator are 128 consecutive
// columns of the output (weight columns, output features), its columns are output rows.  A warp that reads a
// column of the accumulator therefore holds 32 neighbours of one output row and stores them in
// one access, with no transposition on the way out, and the side that varies (tokens of a small batch, rows
// of a weight) takes the accumulator's columns, where tiles of any multiple of 32 are cheap.
#include <algorithm>
#include <atomic>

#include <cudaTypedefs.h>

#include "mx_common.cuh"
#include "tc05.cuh"

namespace rt {

int mx_check_shape(int64_t rows, int64_t cols);
int mx_check_codes(const void* codes, const void* scales);

__device__ unsigned int g_wait_faults;   // waits that ran out; see rt_mx_wait_faults

constexpr int kSms = 148;                 // of a B200; how many clusters run at once is asked of the device
constexpr int kFirstWorker = 4;          // warp 0: loads, 1: products, 2: tensor memory, 3: scales, from 4: conversion and output
constexpr int kConvGroups = 2;           // of four warps each, in the weight gradient's kernel
constexpr int kWgradThreads = 32 * (kFirstWorker + 4 * kConvGroups);
constexpr int kFp4Threads = 32 * (kFirstWorker + 8);
constexpr int kPairGroups = 2;           // of four output warps each
constexpr int kPairThreads = 32 * (kFirstWorker + 4 * kPairGroups);

struct OutMatrix {
  void* p;
  int64_t ld;
  int rows, cols;                        // the accumulator's columns / lanes
  int dtype, accumulate;
  int wide;                              // rows start on 16-byte boundaries
};

template <int D>
__device__ __forceinline__ void put_one(const OutMatrix& o, int64_t at, float v) {
  elem_t<D>* p = static_cast<elem_t<D>*>(o.p) + at;
  *p = of_f32<D>(o.accumulate ? to_f32<D>(*p) + v : v);
}
__device__ __forceinline__ void put_out(const OutMatrix& o, int64_t at, float v) {
  if (o.dtype == RT_BF16) put_one<RT_BF16>(o, at, v);
  else if (o.dtype == RT_F32) put_one<RT_F32>(o, at, v);
  else put_one<RT_F16>(o, at, v);
}
// What is not formed because a wait ran out reads as NaN, so that no such result passes for one: column `col` of the
// output in up to 32 rows from `row`, added to or not.
template <typename T>
__device__ __forceinline__ void fill_column(void* p, int64_t ld, int row, int rows, int col, T v) {
  T* q = static_cast<T*>(p) + (int64_t)row * ld + col;
#pragma unroll 1
  for (int j = 0; j < 32 && row + j < rows; ++j) q[j * ld] = v;
}
__device__ __forceinline__ void put_nan(void* p, int64_t ld, int row, int rows, int col, int cols, int dtype) {
  if (col >= cols) return;
  if (dtype == RT_F32) fill_column<uint32_t>(p, ld, row, rows, col, 0x7FC00000u);
  else fill_column<uint16_t>(p, ld, row, rows, col, dtype == RT_BF16 ? 0x7FC0 : 0x7E00);
}
// 16 columns of the accumulator that this warp holds, to 16 output rows
template <int D>
__device__ __forceinline__ void put_columns(const OutMatrix& o, int row, int col, const uint32_t (&acc)[16]) {
  if (col >= o.cols) return;
  elem_t<D>* p = static_cast<elem_t<D>*>(o.p) + (int64_t)row * o.ld + col;
  const int live = min(16, o.rows - row);
  if (o.accumulate) {
    float old[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) old[j] = j < live ? to_f32<D>(p[j * o.ld]) : 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < live) p[j * o.ld] = of_f32<D>(old[j] + __uint_as_float(acc[j]));
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < live) p[j * o.ld] = of_f32<D>(__uint_as_float(acc[j]));
  }
}

// 32 columns of the accumulator, from this warp's quarter of the lanes, as 32 output rows of 32 values:
// through 2 KB of shared memory that the warp has to itself (fp32 in two halves), so that a lane stores 16
// bytes of one row.  The 16 bytes of a 64-byte row are exchanged by the row's bits 1 and 2, so that the
// eight rows that a transposed store writes lie in different banks.  The instructions of this part bound tiles of
// short sums: with a 16-bit store to each value 8 tokens x 4096 x 4096 took 21.5 us, with pairs rounded together and stored
// transposed 18.6; MXFP4 8192 x 11008 x 4096 156 and 143.  Two squares at a time (19.3, 144) and TMA stores from shared memory were no faster.
template <int D>
__device__ __forceinline__ void put_room(const OutMatrix& o, int row, int col, const elem_t<D>* room) {
  constexpr int kLanes = D == RT_F32 ? 8 : 4, kPer = 16 / (int)sizeof(elem_t<D>), kRows = 32 / kLanes;   // lanes to a row, values to a lane, rows to a store
  const int lane = threadIdx.x & 31, c = col + lane % kLanes * kPer;
  if (row + 4 * kRows <= o.rows && col + 32 <= o.cols) {
    elem_t<D>* p = static_cast<elem_t<D>*>(o.p) + (int64_t)(row + lane / kLanes) * o.ld + c;
    const int64_t hop = kRows * o.ld;
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * kRows + lane / kLanes;
      v[i] = *reinterpret_cast<const uint4*>(room + r * 32 + (D == RT_F32 ? lane % kLanes : lane % kLanes ^ (r >> 1 & 3)) * kPer);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(p + i * hop) = v[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * kRows + lane / kLanes;
    if (row + r < o.rows && c < o.cols) {
      const int chunk = D == RT_F32 ? lane % kLanes : lane % kLanes ^ (r >> 1 & 3);
      const uint4 v = *reinterpret_cast<const uint4*>(room + r * 32 + chunk * kPer);
      elem_t<D>* p = static_cast<elem_t<D>*>(o.p) + (int64_t)(row + r) * o.ld + c;
      if (c + kPer <= o.cols) *reinterpret_cast<uint4*>(p) = v;
      else {
        const elem_t<D>* e = reinterpret_cast<const elem_t<D>*>(&v);
#pragma unroll
        for (int k = 0; k < kPer; ++k)
          if (c + k < o.cols) p[k] = e[k];
      }
    }
  }
}
template <int D>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (D == RT_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <int D>
__device__ __forceinline__ void put_square(const OutMatrix& o, uint32_t tmem, int row, int col, elem_t<D>* room) {
  const int lane = threadIdx.x & 31;
  uint32_t acc[2][16];
  if constexpr (D == RT_F32) {
    tmem_load16(tmem, acc[0]);
    tmem_load16(tmem + 16, acc[1]);
    tmem_wait(acc[0]);
    tmem_wait(acc[1]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < 16; ++j) room[j * 32 + lane] = __uint_as_float(acc[h][j]);
      __syncwarp();
      put_room<D>(o, row + 16 * h, col, room);
      __syncwarp();
    }
  } else {
    tmem_load_fragments(tmem, acc[0]);
    tmem_load_fragments(tmem + (16u << 16), acc[1]);
    tmem_wait(acc[0]);
    tmem_wait(acc[1]);
    const uint32_t to = smem_u32(room) + (lane & 7) * 64 + (((lane >> 3) ^ (lane >> 1 & 3)) << 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {            // eight columns, 32 lanes: four matrices
      uint32_t w[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const uint32_t* p = acc[m >> 1] + 4 * i + 2 * (m & 1);
        w[m] = pack2<D>(__uint_as_float(p[0]), __uint_as_float(p[1]));
      }
      store_transposed(to + i * 512, w[0], w[1], w[2], w[3]);
    }
    __syncwarp();
    put_room<D>(o, row, col, room);
    __syncwarp();
  }
}

// The same added to what the output holds: the sums stay fp32 until they are added, 16 rows at a time.
// What is held is asked for before anything else.  512 tokens x 4096 x 4096, bf16: 34.5 us, value by value from
// the registers 43 (without adding 24); the tile fetched into L2 during the sum made no difference.
template <int D>
__device__ __forceinline__ void add_square(const OutMatrix& o, uint32_t tmem, int row, int col, float* room) {
  constexpr int kPer = 16 / (int)sizeof(elem_t<D>), kLanes = 32 / kPer, kRows = 32 / kLanes, kHops = 16 / kRows;
  const int lane = threadIdx.x & 31, r0 = lane / kLanes, c0 = lane % kLanes * kPer, c = col + c0;
  elem_t<D>* p = static_cast<elem_t<D>*>(o.p) + (int64_t)(row + r0) * o.ld + c;
  const bool full = c + kPer <= o.cols;
  uint4 held[2 * kHops];
#pragma unroll
  for (int i = 0; i < 2 * kHops; ++i)
    held[i] = full && row + i * kRows + r0 < o.rows ? *reinterpret_cast<const uint4*>(p + i * kRows * o.ld) : make_uint4(0, 0, 0, 0);
  uint32_t acc[2][16];
  tmem_load16(tmem, acc[0]);
  tmem_load16(tmem + 16, acc[1]);
  tmem_wait(acc[0]);
  tmem_wait(acc[1]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int j = 0; j < 16; ++j) room[j * 32 + lane] = __uint_as_float(acc[h][j]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kHops; ++i) {
      const int g = h * kHops + i;
      if (row + g * kRows + r0 >= o.rows || c >= o.cols) continue;
      float v[kPer];
#pragma unroll
      for (int k = 0; k < kPer; k += 4) {
        const float4 f = *reinterpret_cast<const float4*>(room + (i * kRows + r0) * 32 + c0 + k);
        v[k] = f.x; v[k + 1] = f.y; v[k + 2] = f.z; v[k + 3] = f.w;
      }
      if (full) {
        const elem_t<D>* e = reinterpret_cast<const elem_t<D>*>(&held[g]);
#pragma unroll
        for (int k = 0; k < kPer; ++k) v[k] += to_f32<D>(e[k]);
        uint4 w;
        if constexpr (D == RT_F32) w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        else w = make_uint4(pack2<D>(v[0], v[1]), pack2<D>(v[2], v[3]), pack2<D>(v[4], v[5]), pack2<D>(v[6], v[7]));
        *reinterpret_cast<uint4*>(p + g * kRows * o.ld) = w;
      } else {
#pragma unroll
        for (int k = 0; k < kPer; ++k)
          if (c + k < o.cols) put_one<D>(o, (int64_t)(row + g * kRows + r0) * o.ld + c + k, v[k]);
      }
    }
    __syncwarp();
  }
}

// The worker warps' part after the last product.  One CTA per tile: straight from tensor memory.
// A cluster per tile (the sum is split over its CTAs): every CTA leaves its part in shared memory, then adds
// up a share of the tile's columns over all of them, always in the order of their ranks.
// `first`, `step`: the cluster's ranks that share this tile.
template <int BN, int WORKERS, bool ADDS>
__device__ __forceinline__ void finish_tile(const OutMatrix& o, uint32_t tmem, int row0, int col0, int splits, int first, int step, float* parts, bool ok) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = warp & 3;
  const bool worker = warp >= kFirstWorker;
  if (worker) {
    constexpr int kGroups = WORKERS / 4;
    const int group = (warp - kFirstWorker) / 4;
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
    if (ok) {
#pragma unroll 1
      for (int c = group * 32; c < BN; c += kGroups * 32) {       // the groups of four warps take 32 columns in turn
        if (splits == 1) {
          if (row0 + c >= o.rows) break;
          if (o.wide && !o.accumulate) {
            float* room = parts + (warp - kFirstWorker) * 512;
            if (o.dtype == RT_BF16) put_square<RT_BF16>(o, lanes + c, row0 + c, col0 + q * 32, reinterpret_cast<uint16_t*>(room));
            else if (o.dtype == RT_F32) put_square<RT_F32>(o, lanes + c, row0 + c, col0 + q * 32, room);
            else put_square<RT_F16>(o, lanes + c, row0 + c, col0 + q * 32, reinterpret_cast<uint16_t*>(room));
            continue;
          }
          if constexpr (ADDS) {
            if (o.wide) {
              float* room = parts + (warp - kFirstWorker) * 512;
              if (o.dtype == RT_BF16) add_square<RT_BF16>(o, lanes + c, row0 + c, col0 + q * 32, room);
              else if (o.dtype == RT_F32) add_square<RT_F32>(o, lanes + c, row0 + c, col0 + q * 32, room);
              else add_square<RT_F16>(o, lanes + c, row0 + c, col0 + q * 32, room);
              continue;
            }
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t acc[16];
          tmem_load16(lanes + c + 16 * h, acc);
          tmem_wait(acc);
          if (splits == 1) {
            if (o.dtype == RT_BF16) put_columns<RT_BF16>(o, row0 + c + 16 * h, col0 + q * 32 + lane, acc);
            else if (o.dtype == RT_F32) put_columns<RT_F32>(o, row0 + c + 16 * h, col0 + q * 32 + lane, acc);
            else put_columns<RT_F16>(o, row0 + c + 16 * h, col0 + q * 32 + lane, acc);
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) parts[(c + 16 * h + j) * 128 + q * 32 + lane] = __uint_as_float(acc[j]);
          }
        }
      }
    } else {
#pragma unroll 1
      for (int c = group * 32; c < BN; c += kGroups * 32) {
        if (splits == 1) put_nan(o.p, o.ld, row0 + c, o.rows, col0 + q * 32 + lane, o.cols, o.dtype);
        else
#pragma unroll 1
          for (int j = 0; j < 32; ++j) parts[(c + j) * 128 + q * 32 + lane] = __uint_as_float(0x7FC00000u);
      }
    }
    tc_fence_before();
  }
  if (splits > 1) {
    __syncwarp();
    cluster_sync();
    if (worker) {
      const int rank = ((int)cluster_rank() - first) / step;
      const uint32_t base = smem_u32(parts);
      for (int e = threadIdx.x - kFirstWorker * 32; e < (BN + splits - 1) / splits * 32; e += WORKERS * 32) {   // four lanes of one column
        const int c = rank + (e >> 5) * splits, f = (e & 31) * 4, col = col0 + f;
        if (c >= BN) break;
        float4 v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r < splits) v[r] = load_peer(base + (uint32_t)(c * 128 + f) * 4, first + r * step);
        float sum[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
        for (int r = 1; r < 8; ++r)
          if (r < splits) { sum[0] += v[r].x; sum[1] += v[r].y; sum[2] += v[r].z; sum[3] += v[r].w; }
        if (row0 + c < o.rows)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (col + j < o.cols) put_out(o, (int64_t)(row0 + c) * o.ld + col + j, sum[j]);
      }
    }
    __syncwarp();
    cluster_sync();
  }
}

// ------------------------------------------------------------------------------- weight gradient
// D[k, n] = sum over tokens of value(k, t) * grad(t, n).  Both operands lie with the token as the
// slow index, so both are MN-major; a step takes 64 tokens.  The gradient's tile comes by TMA
// ready for the tensor core; the codes' tile (8 KB) comes by TMA as bytes, the worker warps turn
// it into bf16 (exact: a code times a power of two) in the swizzled layout.  fp32 and fp16
// gradients arrive as up to three bf16 pieces that add up to them; the pieces are further steps of the same sum.
//
// PAIR: two CTAs (ranks 2j and 2j + 1 of a cluster) make one tile of 256 features x BN, each with its own
// 128 features and half of the gradient's columns, so that the gradient's tile is fetched and read half as
// often: one CTA's 40 KB a step at 128 x 256 keep the L2 busier than the tensor core.  Rank 2j issues the
// products; both CTAs' workers arrive at its barrier.
//
// What bounds it: at BN = 512 (all of tensor memory; a step's converted tile serves two products) the
// tensor core, 472-482 us at 8192 x 4096 x 11008 = 1530-1560 TFLOP/s (taking out the conversion changed nothing); below that
// the conversion, some 0.4 us a step (8192 codes; four integer operations to a pair, and the pipe
// takes a warp in two clocks): 18.8 us at 2048 x 1024 x 4096, 14.8 at 16384 x 256 x 512.
// The sums are what the tensor core makes of them: it cuts the bits that do not fit, so that an fp32 result comes out
// a little small.  Off by (relative norm, normal data, 4096 x 4096 outputs) 2e-7 at 1024 tokens, 2.7e-6 at 8192, 7e-6 at 16384, as
// the library's bf16 product with fp32 results is to the digit; where the sum is split, as the shorter sums are.
constexpr int kTok = 64;

template <int BN, bool PAIR>
struct WgradSmem {
  static constexpr int kCols = PAIR ? BN / 2 : BN;                // gradient columns that this CTA fetches
  static constexpr int kCodes = 128 * kTok, kA = 128 * kTok * 2, kB = kCols * kTok * 2, kScales = kTok * 4;
  static constexpr int kStage = kCodes + kA + kB + kScales;
  static constexpr int kStages = kCols == 256 ? 4 : kCols == 128 ? 5 : 6;
  static constexpr int kBytes = kStages * kStage + 1024 + 256;   // alignment, barriers
  static constexpr int kN = BN > 256 ? 256 : BN;                  // columns to a product; BN / kN products share A
};

struct WgradArgs {
  const uint8_t* scales;
  int64_t ld_scales;
  int tokens;
  int token_steps, pieces, splits;
  int k_tiles, n_tiles;                   // k_tiles: of 256 features with PAIR, else of 128
  int64_t part;                           // 0, or bytes between the parts of a sum that another kernel joins (see join_parts_kernel)
  OutMatrix out;
};

// Two codes in the low bytes of the halves of a word -> two bf16 numbers code * 2^(byte - 133).  With
// code = low7 - 128 * (top bit), (128 + low7) * 2^m and (128 + 128 * (top bit)) * 2^m are bf16 numbers made by
// setting and adding bits to k = the bits of 128 * 2^m, m = byte - 133, and their difference is exact.  k is
// (byte + 1) << 7, which has an exponent for every byte up to 252; a warp that meets a larger one
// (values from 2^119 on, or NaN) multiplies by the scale instead.
__device__ __forceinline__ uint32_t bf16x2_of_codes(uint32_t w, uint32_t k) {
  const uint32_t x = (w & 0x007F007Fu) | k, y = (w & 0x00800080u) + k;
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
  return *reinterpret_cast<const uint32_t*>(&v);
}
constexpr uint32_t kByteOfOne = 133;     // the scale byte of 2^0
__device__ __forceinline__ uint32_t scaled(uint32_t v, uint32_t byte) {
  const uint32_t h = byte == 255u ? 0x7FC0u : byte >= 7u ? (byte - 6u) << 7 : 1u << byte, w = h | h << 16;   // 2^(byte - 133)
  const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&w));
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <int BN, bool PAIR>
__global__ void __launch_bounds__(kWgradThreads, 1)
mx_weight_grad_kernel(const __grid_constant__ CUtensorMap map_codes, const __grid_constant__ CUtensorMap map_grad, const WgradArgs a) {
  using S = WgradSmem<BN, PAIR>;
  static_assert(BN > 256 || BN * 512 <= S::kStages * S::kStage, "a part of a split tile");
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t tile_a = base, tile_b = tile_a + S::kStages * S::kA, codes = tile_b + S::kStages * S::kB;
  const uint32_t scales = codes + S::kStages * S::kCodes, bars = scales + S::kStages * S::kScales;
  const uint32_t full = bars, empty = bars + 8 * S::kStages, conv = empty + 8 * S::kStages, done = conv + 8 * S::kStages, slot = done + 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // tiles: groups of eight along n, k inside: the CTAs that run together share few tiles of either side
  constexpr int kCtas = PAIR ? 2 : 1;
  const int in_cluster = blockIdx.x % (a.splits * kCtas), side = PAIR ? in_cluster & 1 : 0, split = in_cluster / kCtas;
  const int tile = blockIdx.x / (a.splits * kCtas);
  const int per_group = 8 * a.k_tiles, group = tile / per_group, width = min(8, a.n_tiles - 8 * group);
  const int in_group = tile - group * per_group;
  const int n0 = (group * 8 + in_group % width) * BN, k0 = (in_group / width * kCtas + side) * 128;
  const int64_t steps = (int64_t)a.token_steps * a.pieces;
  const int first = (int)(steps * split / a.splits), count = (int)(steps * (split + 1) / a.splits) - first;
  const uint32_t leader = PAIR ? cluster_rank() & ~1u : 0u;

  if (warp == 0 && elect_one()) {
    prefetch_map(&map_codes);
    prefetch_map(&map_grad);
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(full + 8 * s, 1 + 32);       // the loads, and warp 3's lanes
      mbar_init(empty + 8 * s, 1 + 4 * (kConvGroups - 1));      // the products, and the warps that have only looked at the step
      mbar_init(conv + 8 * s, 4 * kCtas);    // the four warps of a step, of both CTAs
    }
    mbar_init(done, 1);
    fence_barrier_init();
  }
  constexpr int kColumns = BN, kHalfN = S::kN / kCtas;     // columns of one product that this CTA holds
  if (warp == 2) tmem_alloc<PAIR>(slot, kColumns);
  __syncthreads();
  if constexpr (PAIR) cluster_sync();        // the other CTA's barriers are there
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + (slot - base));
  bool ok = true;

  if (warp == 0) {
    if (elect_one()) {
      int piece = first / a.token_steps, t = first % a.token_steps, i = 0;
      for (; i < count; ++i) {
        const int s = i % S::kStages;
        if (!(ok = mbar_wait(empty + 8 * s, ((i / S::kStages) & 1) ^ 1))) break;
        mbar_expect(full + 8 * s, S::kCodes + S::kB);
        tma_load_2d(&map_codes, codes + s * S::kCodes, full + 8 * s, k0, t * kTok);
#pragma unroll
        for (int j = 0; j < S::kCols / 64; ++j)
          tma_load_3d(&map_grad, tile_b + s * S::kB + j * 8192, full + 8 * s, n0 + (j * 64 / kHalfN) * S::kN + side * kHalfN + j * 64 % kHalfN, t * kTok, piece);
        if (++t == a.token_steps) { t = 0; ++piece; }
      }
      if (!ok)   // the loads in flight still write to this CTA's memory
        for (int j = 0; j < S::kStages && j < i; ++j) {
          const int latest = i - 1 - (i - 1 - j) % S::kStages;       // the last step that used stage j
          mbar_wait(full + 8 * j, (latest / S::kStages) & 1);
        }
    }
  } else if (warp == 1) {
    if (side == 0 && elect_one()) {
      constexpr uint32_t idesc = idesc_bf16_mn(128 * kCtas, S::kN);
      const uint16_t both = (uint16_t)(3u << leader);
      for (int i = 0; i < count; ++i) {
        const int s = i % S::kStages, phase = (i / S::kStages) & 1;
        if (!(ok = mbar_wait(full + 8 * s, phase) && mbar_wait(conv + 8 * s, phase))) break;
        tc_fence_after();
        const uint64_t da = tile_desc(tile_a + s * S::kA, 8192, 1024), db = tile_desc(tile_b + s * S::kB, 8192, 1024);
#pragma unroll
        for (int kk = 0; kk < kTok / 16; ++kk)
#pragma unroll
          for (int j = 0; j < BN / S::kN; ++j)
            mma_bf16<PAIR>(tmem + j * S::kN, da + kk * (2048 >> 4), db + ((j * kHalfN * kTok * 2 + kk * 2048) >> 4), idesc, i > 0 || kk > 0);
        tc_commit<PAIR>(empty + 8 * s, both);
      }
      if (ok) tc_commit<PAIR>(done, both);   // otherwise the workers' wait runs out too, and they leave NaN
    }
  } else if (warp == 3) {
    // the scales of a step: one word (four blocks) to a token
    const uint8_t* sc = a.scales + (k0 >> 5);
    const bool some = (k0 >> 5) < a.ld_scales;      // the second CTA of the last pair may have nothing
    int t = first % a.token_steps;
    for (int i = 0; i < count; ++i) {
      const int s = i % S::kStages;
      if (!(ok = mbar_wait_warp(empty + 8 * s, ((i / S::kStages) & 1) ^ 1))) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int token = t * kTok + h * 32 + lane;
        const bool live = some && token < a.tokens;
        copy4(scales + s * S::kScales + (h * 32 + lane) * 4, live ? sc + token * a.ld_scales : a.scales, live);
      }
      copies_arrive(full + 8 * s);
      if (++t == a.token_steps) t = 0;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp >= kFirstWorker) {
    // Two groups of four warps take the steps in turn (four groups were no faster); 64 codes to a thread, 16 of them (a chunk of the
    // codes, two of the bf16 tile) at a time.  Lanes 0-3 and 4-7, and so on, have tokens that differ in bits 0 and 2: with
    // both tiles' chunks exchanged by the token's low bits (128-byte swizzle), eight lanes then read eight
    // different chunks of a row and write eight different ones.
    const int w = warp & 3, sub = lane & 3, pair = lane >> 3, low = lane & 4 ? pair ^ 5 : pair;      // low: token & 7
    const int mine = (warp - kFirstWorker) >> 2;
    for (int i = 0; i < count; ++i) {
      const int s = i % S::kStages, phase = (i / S::kStages) & 1;
      // Every phase in turn: one that was left out could be taken for the next but one.  The group whose step it is
      // not says that it has seen the phase: the stage is not filled anew before, so none can pass unseen.  (Said to the products
      // instead, over the pair, it took 10 ns a step more.)
      if (!(ok = mbar_wait_warp(full + 8 * s, phase))) break;
      if (i % kConvGroups != mine) {
        if (lane == 0) mbar_arrive(empty + 8 * s);
        continue;
      }
      const uint8_t* in = smem + (codes - base) + s * S::kCodes + (w * 16 + low) * 128;
      const uint8_t* sc = smem + (scales - base) + s * S::kScales + (w * 16 + low) * 4;
      uint8_t* out = smem + (tile_a - base) + s * S::kA + (w * 16 + low) * 128;
      uint4 c[4];
      uint32_t byte[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) {      // token groups h / 2, feature halves h % 2
        c[h] = *reinterpret_cast<const uint4*>(in + (h >> 1) * 1024 + ((((h & 1) * 4 + sub) ^ low) << 4));
        byte[h] = sc[(h >> 1) * 32 + (h & 1) * 2 + (sub >> 1)];
      }
      const bool slow = __any_sync(0xFFFFFFFFu, max(max(byte[0], byte[1]), max(byte[2], byte[3])) > 252u);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const uint32_t k = ((slow ? kByteOfOne : byte[h]) + 1u) * 0x00800080u;
        const uint32_t u[4] = {c[h].x, c[h].y, c[h].z, c[h].w};
        uint32_t v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[2 * j] = bf16x2_of_codes(__byte_perm(u[j], 0u, 0x4140), k);
          v[2 * j + 1] = bf16x2_of_codes(__byte_perm(u[j], 0u, 0x4342), k);
        }
        if (slow) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = scaled(v[j], byte[h]);
        }
        uint8_t* row = out + (h >> 1) * 1024 + (h & 1) * 8192;
        *reinterpret_cast<uint4*>(row + (((sub * 2) ^ low) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<uint4*>(row + (((sub * 2 + 1) ^ low) << 4)) = make_uint4(v[4], v[5], v[6], v[7]);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) mbar_arrive_at(conv + 8 * s, leader);
        else mbar_arrive(conv + 8 * s);
      }
    }
    ok = mbar_wait_warp(done, 0) && ok;
    tc_fence_after();
  }
  __syncwarp();
  if (!ok) atomicAdd(&g_wait_faults, 1u);
  OutMatrix o = a.out;
  if (a.part) o.p = static_cast<uint8_t*>(o.p) + split * a.part;
  finish_tile<BN, 4 * kConvGroups, true>(o, tmem, n0, k0, a.part ? 1 : a.splits, side, kCtas, reinterpret_cast<float*>(smem), ok);
  __syncthreads();
  if constexpr (PAIR) cluster_meet();        // the pair's products read both CTAs' memory, its barriers are in both
  if (warp == 2) tmem_free<PAIR>(tmem, kColumns);
}

// Few tiles and a long sum: more splits than a cluster has CTAs, each leaving its part of the output in
// fp32, and this kernel adds them up in their order.  Four columns to a thread.  65536 x 256 x 512: 25 us
// (in clusters of eight, which run 15 at a time, 54), 16384 x 256 x 512: 14.8 (18).  18 parts of 256 x 512 take it 3 us, bound by
// the latency of its loads.
__global__ void __launch_bounds__(256)
join_parts_kernel(const float4* __restrict__ parts, const int64_t quads, const int splits, const FastDiv per_row, const OutMatrix o) {
  const uint32_t q = blockIdx.x * 256 + threadIdx.x;
  if (q >= quads) return;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int s = 0; s < splits; ++s) {
    const float4 v = __ldcs(parts + s * quads + q);
    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
  }
  uint32_t r, c;
  per_row.split(q, r, c);
  const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if ((int)c * 4 + j < o.cols) put_out(o, (int64_t)r * o.ld + c * 4 + j, v[j]);
}

// A gradient that the tensor maps cannot take as it is (fp32, fp16, rows that do not start on 16-byte
// boundaries) as bf16 planes whose sum it is (down to 2^-133, the last place of a bf16 number): the
// leading 8 bits of each value's mantissa, the next 8, the rest.  Cut, not rounded, so that nothing overflows; an infinity or a NaN is in the first plane alone.
// 4096 x 4096 fp32: 24 us, bound by the integer pipe (66 %) and memory (67 MB read, 100 written); the planes cost more in what follows, the
// codes being widened once for each: 4096 x 4096 x 1024 takes 103-115 us from fp32, 78-82 from fp16.
// Eight values of a row to a thread, of two rows, planes of np = n rounded up to eight columns.
template <int D, int P, bool VEC>
__global__ void __launch_bounds__(256)
spread_gradient_kernel(const Matrix g, const FastDiv upr, const int64_t tokens, const int n, uint16_t* __restrict__ planes) {
  uint32_t group, c8;
  upr.split(blockIdx.x * 256 + threadIdx.x, group, c8);
  const int64_t row = (int64_t)group * 2, total = tokens * upr.d * 8;
  Raw8<D> raw[2];
  load_rows<D, VEC>(g, row, 1, (int)c8 * 8, n, tokens, raw);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (row + r >= tokens) break;
    uint16_t* out = planes + (row + r) * upr.d * 8 + c8 * 8;
    if constexpr (P == 1) {
      *reinterpret_cast<uint4*>(out) = raw[r].w[0];
    } else {
      float v[8];
      unpack<D>(raw[r], v);
      uint32_t b[8];
      bool odd[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        b[k] = __float_as_uint(v[k]);
        odd[k] = (b[k] & 0x7F800000u) == 0x7F800000u;
        if (odd[k] && (b[k] & 0x7FFFFFu)) b[k] = 0x7FC00000u;
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        *reinterpret_cast<uint4*>(out + p * total) = make_uint4(__byte_perm(b[0], b[1], 0x7632), __byte_perm(b[2], b[3], 0x7632),
                                                                __byte_perm(b[4], b[5], 0x7632), __byte_perm(b[6], b[7], 0x7632));
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          v[k] = odd[k] ? 0.f : v[k] - __uint_as_float(b[k] & 0xFFFF0000u);
          b[k] = __float_as_uint(v[k]);
        }
      }
    }
  }
}
template <int D, int P>
static void run_spread(const void* g, int64_t ld, int64_t tokens, int64_t n, void* planes, cudaStream_t st) {
  const FastDiv upr = FastDiv::of((uint32_t)((n + 7) / 8));
  const unsigned nb = (unsigned)(((uint64_t)((tokens + 1) / 2) * upr.d + 255) / 256);
  auto k = aligned16(g, ld, (int)sizeof(elem_t<D>)) ? spread_gradient_kernel<D, P, true> : spread_gradient_kernel<D, P, false>;
  k<<<nb, 256, 0, st>>>({g, ld}, upr, tokens, (int)n, (uint16_t*)planes);
}

// ---------------------------------------------------------------------------------- fp4 product
// D[n, m] = sum over k of b[n, k] * a[m, k]: the 128 lanes are rows of b (output features), the
// columns rows of a (tokens).  Codes go from global memory to the tensor core as they are stored: a
// step is 256 columns, 128 bytes of a row, K-major.  The scales lie in global memory in the order
// that tensor memory wants, so a row tile's scales of a step are one bulk copy to shared memory and
// two copies (one per 128 columns) to tensor memory, where each stage has columns of its own.
// The product takes a tile's scales from where a scale tile begins (an odd column of tensor memory
// is a misaligned address to it), so narrow tiles serve only matrices of a single tile of rows.
// One token against 11008 x 4096: 8.2-8.6 us (24 MB at 2.8-2.9 TB/s).  What bounds it there is the chain of a step, 0.34 us:
// scales, four products that add to the same sums, release; twice the loads under way changed nothing.
constexpr int kStepK = 256;

template <int BN>
struct Fp4Smem {
  static constexpr int kA = 128 * 128, kB = BN * 128, kScale = 1024;
  static constexpr int kStage = kA + kB + 2 * kScale;
  static constexpr int kStages = BN == 128 ? 3 : BN == 64 ? 4 : 5;   // two CTAs to an SM
  static constexpr int kBytes = kStages * kStage + 1024 + 256;
  static constexpr int kColumns = BN + 16 * kStages <= 128 ? 128 : 256;
};

struct Fp4Args {
  const uint8_t* a_scales;
  const uint8_t* b_scales;
  int k_padded, steps, ktiles, splits;
  int n_tiles, m_tiles;
  OutMatrix out;
};

template <int BN>
__global__ void __launch_bounds__(kFp4Threads, 2)
mx_fp4_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Fp4Args a) {
  using S = Fp4Smem<BN>;
  static_assert(BN * 512 <= S::kStages * S::kStage, "a part of a split tile");
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t tile_b = base, tile_a = tile_b + S::kStages * S::kA, scale_b = tile_a + S::kStages * S::kB;   // b's rows are the lanes
  const uint32_t scale_a = scale_b + S::kStages * S::kScale, bars = scale_a + S::kStages * S::kScale;
  const uint32_t full = bars, empty = bars + 8 * S::kStages, done = empty + 8 * S::kStages, slot = done + 8;
  const int warp = threadIdx.x >> 5;

  const int tile = blockIdx.x / a.splits, rank = blockIdx.x % a.splits;
  const int per_group = 8 * a.n_tiles, group = tile / per_group, width = min(8, a.m_tiles - 8 * group);
  const int in_group = tile - group * per_group;
  const int m0 = (group * 8 + in_group % width) * BN, nt = in_group / width, n0 = nt * 128;
  const int first = (int)((int64_t)a.steps * rank / a.splits), last = (int)((int64_t)a.steps * (rank + 1) / a.splits);

  if (warp == 0 && elect_one()) {
    prefetch_map(&map_a);
    prefetch_map(&map_b);
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1);
    }
    mbar_init(done, 1);
    fence_barrier_init();
  }
  if (warp == 2) tmem_alloc<false>(slot, S::kColumns);
  __syncthreads();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + (slot - base));
  bool ok = true;

  if (warp == 0) {
    if (elect_one()) {
      const uint8_t* sb = a.b_scales + (int64_t)nt * a.ktiles * 512;
      const uint8_t* sa = a.a_scales + (int64_t)(m0 >> 7) * a.ktiles * 512;
      int i = 0;
      for (int it = first; it < last; ++it, ++i) {
        const int s = i % S::kStages;
        if (!(ok = mbar_wait(empty + 8 * s, ((i / S::kStages) & 1) ^ 1))) break;
        const uint32_t bytes = 512u * min(2, a.ktiles - 2 * it);
        mbar_expect(full + 8 * s, S::kA + S::kB + 2 * bytes);
        tma_load_2d(&map_b, tile_b + s * S::kA, full + 8 * s, it * 128, n0);
        tma_load_2d(&map_a, tile_a + s * S::kB, full + 8 * s, it * 128, m0);
        bulk_load(scale_b + s * S::kScale, sb + (int64_t)it * 1024, bytes, full + 8 * s);
        bulk_load(scale_a + s * S::kScale, sa + (int64_t)it * 1024, bytes, full + 8 * s);
      }
      if (!ok)   // the loads in flight still write to this CTA's memory
        for (int j = 0; j < S::kStages && j < i; ++j) {
          const int latest = i - 1 - (i - 1 - j) % S::kStages;
          mbar_wait(full + 8 * j, (latest / S::kStages) & 1);
        }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      for (int i = 0; i < last - first; ++i) {
        const int s = i % S::kStages, it = first + i;
        if (!(ok = mbar_wait(full + 8 * s, (i / S::kStages) & 1))) break;
        tc_fence_after();
        const uint32_t sf = tmem + BN + 16 * s;
        const int halves = min(2, a.ktiles - 2 * it), products = min(4, (a.k_padded - it * kStepK + 63) / 64);
        for (int h = 0; h < halves; ++h) {
          copy_scales<false>(sf + 4 * h, plain_desc(scale_b + s * S::kScale + 512 * h, 128, 128));
          copy_scales<false>(sf + 8 + 4 * h, plain_desc(scale_a + s * S::kScale + 512 * h, 128, 128));
        }
        const uint64_t db = tile_desc(tile_b + s * S::kA, 16, 1024), da = tile_desc(tile_a + s * S::kB, 16, 1024);
        for (int kk = 0; kk < products; ++kk)
          mma_mxfp4<false>(tmem, db + kk * 2, da + kk * 2, kk & 1 ? idesc_mxfp4(128, BN, 1) : idesc_mxfp4(128, BN, 0), sf + 4 * (kk >> 1),
                    sf + 8 + 4 * (kk >> 1), i > 0 || kk > 0);
        tc_commit<false>(empty + 8 * s);
      }
      if (ok) tc_commit<false>(done);        // otherwise the workers' wait runs out too, and they leave NaN
    }
  } else if (warp >= kFirstWorker) {
    ok = mbar_wait_warp(done, 0);
    tc_fence_after();
  }
  __syncwarp();
  if (!ok) atomicAdd(&g_wait_faults, 1u);
  finish_tile<BN, 8, false>(a.out, tmem, m0, n0, a.splits, 0, 1, reinterpret_cast<float*>(smem), ok);
  __syncthreads();
  if (warp == 2) tmem_free<false>(tmem, S::kColumns);
}

// Large products: pairs of CTAs stay and take tile after tile, 256 rows of b (128 to a CTA) x 384 rows of a
// (192 to a CTA), as a product of 256 columns and one of 128 per 64 columns of the sum.  What bounds
// the small tiles above is the way from L2: 34 KB per CTA for 256 clocks of products at 128 x 128,
// here 44 KB for 768.  384 columns of sums and four stages of scales (8 columns of b's, 24 of a's) fill
// tensor memory, so a tile's output is not overlapped with the next one's products, but its loads are.
// 8192 x 11008 x 4096: 143 us (5.2 PFLOP/s), 8192 x 8192 x 8192: 188 us (5.8); a step takes 0.5 us, of which the
// products are 0.4, and a tile's start and output 3.
// Every CTA needs the scales of all 384 rows of a.  Both CTAs' loads report to the first one's barrier (told
// by a warp of the second instead, a step took 550 ns); the first issues all copies and products.
struct PairSmem {
  static constexpr int kLanes = 128 * 128, kRows1 = 128 * 128, kRows2 = 64 * 128, kLaneScales = 1024, kRowScales = 3 * 1024;
  static constexpr int kStage = kLanes + kRows1 + kRows2 + kLaneScales + kRowScales;
  static constexpr int kStages = 4, kRoom = 4 * kPairGroups * 2048;
  static constexpr int kBytes = kStages * kStage + kRoom + 1024 + 256;
  static constexpr int kTileRows = 384, kSums = 384, kScaleColumns = 32;
};

__global__ void __launch_bounds__(kPairThreads, 1)
mx_fp4_pair_kernel(const __grid_constant__ CUtensorMap map_a1, const __grid_constant__ CUtensorMap map_a2, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb, const Fp4Args a) {
  using S = PairSmem;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t tile_b = base, tile_a1 = tile_b + S::kStages * S::kLanes, tile_a2 = tile_a1 + S::kStages * S::kRows1;
  const uint32_t scale_b = tile_a2 + S::kStages * S::kRows2, scale_a = scale_b + S::kStages * S::kLaneScales;
  const uint32_t room = scale_a + S::kStages * S::kRowScales, bars = room + S::kRoom;
  const uint32_t full = bars, empty = full + 8 * S::kStages, done = empty + 8 * S::kStages, drained = done + 8, slot = drained + 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, side = blockIdx.x & 1;
  const int tiles = a.n_tiles * a.m_tiles, pairs = gridDim.x >> 1;

  if (warp == 0 && elect_one()) {
    prefetch_map(&map_a1);
    prefetch_map(&map_a2);
    prefetch_map(&map_b);
    prefetch_map(&map_sa);
    prefetch_map(&map_sb);
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(full + 8 * s, 1);            // the first CTA's: expects both CTAs' bytes
      mbar_init(empty + 8 * s, 1);
    }
    mbar_init(done, 1);
    mbar_init(drained, 2 * 4 * kPairGroups); // the output warps of both CTAs
    fence_barrier_init();
  }
  if (warp == 2) tmem_alloc<true>(slot, 512);
  __syncthreads();
  cluster_sync();                            // the other CTA's barriers are there
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + (slot - base));
  bool ok = true;

  // tile t: eight tiles of a's rows side by side, b's inside
  auto place = [&](int t, int& m0, int& n0) {
    const int per_group = 8 * a.n_tiles, group = t / per_group, width = min(8, a.m_tiles - 8 * group), in = t - group * per_group;
    m0 = (group * 8 + in % width) * S::kTileRows;
    n0 = in / width * 256;
  };

  if (warp == 0) {
    if (elect_one()) {
      int i = 0;                             // steps so far, over all tiles
      for (int t = blockIdx.x >> 1; t < tiles && ok; t += pairs) {
        int m0, n0;
        place(t, m0, n0);
        const int row = n0 + side * 128;
        for (int k = 0; k < a.steps; ++k, ++i) {
          const int s = i % S::kStages;
          if (!(ok = mbar_wait(empty + 8 * s, ((i / S::kStages) & 1) ^ 1))) break;
          if (side == 0) mbar_expect(full + 8 * s, 2 * S::kStage);
          const uint32_t bar = address_at(full + 8 * s, 0);
          tma_load_2d_pair(&map_b, tile_b + s * S::kLanes, bar, k * 128, row);
          tma_load_2d_pair(&map_a1, tile_a1 + s * S::kRows1, bar, k * 128, m0 + side * 128);
          tma_load_2d_pair(&map_a2, tile_a2 + s * S::kRows2, bar, k * 128, m0 + 256 + side * 64);
          tma_load_2d_pair(&map_sb, scale_b + s * S::kLaneScales, bar, k * 256, row >> 7);
          tma_load_2d_pair(&map_sa, scale_a + s * S::kRowScales, bar, k * 256, m0 >> 7);
        }
      }
      // If a wait ran out, loads may still be on their way to both CTAs' memory; all of them report to the first CTA's
      // barriers, which it waits for (again with the limit) before the pair's last barrier lets either end.
      if (!ok && side == 0)
        for (int j = 0; j < S::kStages && j < i; ++j) {
          const int latest = i - 1 - (i - 1 - j) % S::kStages;
          mbar_wait(full + 8 * j, (latest / S::kStages) & 1);
        }
    }
  } else if (warp == 1) {
    if (side == 0 && elect_one()) {
      int i = 0, n = 0;
      for (int t = blockIdx.x >> 1; t < tiles && ok; t += pairs, ++n) {
        if (n > 0 && !(ok = mbar_wait(drained, (n - 1) & 1))) break;
        for (int k = 0; k < a.steps; ++k, ++i) {
          const int s = i % S::kStages;
          if (!(ok = mbar_wait(full + 8 * s, (i / S::kStages) & 1))) break;
          tc_fence_after();
          const uint32_t sf = tmem + S::kSums + S::kScaleColumns * s;
          const int halves = min(2, a.ktiles - 2 * k), products = min(4, (a.k_padded - k * kStepK + 63) / 64);
          for (int h = 0; h < halves; ++h) {
            copy_scales<true>(sf + 4 * h, plain_desc(scale_b + s * S::kLaneScales + 512 * h, 128, 128));
#pragma unroll
            for (int r = 0; r < 3; ++r)
              copy_scales<true>(sf + 8 + 12 * h + 4 * r, plain_desc(scale_a + s * S::kRowScales + 1024 * r + 512 * h, 128, 128));
          }
          const uint64_t db = tile_desc(tile_b + s * S::kLanes, 16, 1024), d1 = tile_desc(tile_a1 + s * S::kRows1, 16, 1024), d2 = tile_desc(tile_a2 + s * S::kRows2, 16, 1024);
          for (int kk = 0; kk < products; ++kk) {
            const uint32_t sb = sf + 4 * (kk >> 1), sa = sf + 8 + 12 * (kk >> 1);
            mma_mxfp4<true>(tmem, db + kk * 2, d1 + kk * 2, kk & 1 ? idesc_mxfp4(256, 256, 1) : idesc_mxfp4(256, 256, 0), sb, sa, k > 0 || kk > 0);
            mma_mxfp4<true>(tmem + 256, db + kk * 2, d2 + kk * 2, kk & 1 ? idesc_mxfp4(256, 128, 1) : idesc_mxfp4(256, 128, 0), sb, sa + 8, k > 0 || kk > 0);
          }
          tc_commit<true>(empty + 8 * s, 3);
        }
        if (ok) tc_commit<true>(done, 3);    // otherwise the workers' wait runs out too, and they leave NaN from this tile on
      }
    }
  } else if (warp >= kFirstWorker) {
    const int q = warp & 3, group = (warp - kFirstWorker) >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
    float* space = reinterpret_cast<float*>(smem + (room - base)) + (warp - kFirstWorker) * 512;
    int n = 0;
    for (int t = blockIdx.x >> 1; t < tiles; t += pairs, ++n) {
      int m0, n0;
      place(t, m0, n0);
      const int col = n0 + side * 128 + q * 32;
      if (!(ok = ok && mbar_wait_warp(done, n & 1))) {
#pragma unroll 1
        for (int c = group * 32; c < S::kTileRows; c += 32 * kPairGroups) put_nan(a.out.p, a.out.ld, m0 + c, a.out.rows, col + lane, a.out.cols, a.out.dtype);
        continue;
      }
      tc_fence_after();
#pragma unroll 1
      for (int c = group * 32; c < S::kTileRows && m0 + c < a.out.rows; c += 32 * kPairGroups) {
        if (a.out.wide) {
          if (a.out.dtype == RT_BF16) put_square<RT_BF16>(a.out, lanes + c, m0 + c, col, reinterpret_cast<uint16_t*>(space));
          else if (a.out.dtype == RT_F32) put_square<RT_F32>(a.out, lanes + c, m0 + c, col, space);
          else put_square<RT_F16>(a.out, lanes + c, m0 + c, col, reinterpret_cast<uint16_t*>(space));
          continue;
        }
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          uint32_t acc[16];
          tmem_load16(lanes + c + 16 * h, acc);
          tmem_wait(acc);
          if (a.out.dtype == RT_BF16) put_columns<RT_BF16>(a.out, m0 + c + 16 * h, col + lane, acc);
          else if (a.out.dtype == RT_F32) put_columns<RT_F32>(a.out, m0 + c + 16 * h, col + lane, acc);
          else put_columns<RT_F16>(a.out, m0 + c + 16 * h, col + lane, acc);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_at(drained, 0);
    }
  }
  __syncwarp();
  if (!ok) atomicAdd(&g_wait_faults, 1u);
  tc_fence_before();
  __syncthreads();
  cluster_sync();                            // the products read both CTAs' memory, the barriers are in both
  if (warp == 2) tmem_free<true>(tmem, 512);
}

static int check_out(const void* out, int dtype, int64_t cols, int64_t ld) {
  if (!out) return fail(RT_E_NULL, "out must be non-null");
  if (!dtype_ok(dtype)) return fail(RT_E_DTYPE, "dtype code must be 0 (bf16), 1 (f32) or 2 (f16)");
  if (ld < cols || ld > ((int64_t)1 << 40)) return fail(RT_E_SIZE, "row stride of out must be >= cols and at most 2^40");
  if ((uintptr_t)out % dtype_size(dtype)) return fail(RT_E_ALIGN, "out is not aligned to its element size");
  return 0;
}
static int launched() {
  stats().kernel_launches.fetch_add(1, std::memory_order_relaxed);
  RT_CUDA(cudaGetLastError());
  return 0;
}


static PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
  static std::atomic<void*> fn{nullptr};
  void* p = fn.load(std::memory_order_acquire);
  if (!p) {
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
      return nullptr;
    fn.store(p, std::memory_order_release);
  }
  return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
}
// dims and box from the innermost dimension; strides (bytes) of all but the innermost
static int make_map(CUtensorMap* map, CUtensorMapDataType type, const void* p, int rank, const uint64_t* dims, const uint64_t* strides,
                    const uint32_t* box, CUtensorMapSwizzle swizzle) {
  auto encode = map_encoder();
  if (!encode) { cudaGetLastError(); return fail(RT_E_DEVICE, "the driver has no cuTensorMapEncodeTiled"); }
  const cuuint32_t ones[3] = {1, 1, 1};
  const auto fill = [&] {
    return encode(map, type, (cuuint32_t)rank, const_cast<void*>(p), reinterpret_cast<const cuuint64_t*>(dims),
                  reinterpret_cast<const cuuint64_t*>(strides), box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = fill();
  if (r == CUDA_ERROR_INVALID_CONTEXT || r == CUDA_ERROR_NOT_INITIALIZED) {   // a thread's first call (autograd's, for one): the runtime has not bound the device's context yet
    int device = 0;
    RT_CUDA(cudaGetDevice(&device));
    RT_CUDA(cudaSetDevice(device));
    r = fill();
  }
  if (r != CUDA_SUCCESS) return fail(RT_E_CONFIG, "cuTensorMapEncodeTiled failed: " + std::to_string((int)r));
  return 0;
}

// Launch a tensor-core kernel as clusters of `cluster` CTAs.  Its shared memory is raised once per
// device and kernel.
template <typename K, typename... Args>
static int launch_tc(K kernel, std::atomic<uint64_t>& raised, int threads, int smem, int64_t ctas, int cluster, cudaStream_t st, Args... args) {
  int device = 0;
  RT_CUDA(cudaGetDevice(&device));
  if (device >= 64 || !(raised.load(std::memory_order_acquire) >> device & 1)) {
    RT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    RT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    if (device < 64) raised.fetch_or(1ull << device, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)cluster;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  RT_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  stats().kernel_launches.fetch_add(1, std::memory_order_relaxed);
  return 0;
}

// How many clusters of `cluster` CTAs of a kernel the device runs at once: fewer than its SMs would
// hold, since a cluster stays within a group of SMs (15 of eight CTAs, 33 of four on 148 SMs).  Asked once
// per device, kernel and size.
template <typename K>
static int clusters_at_once(K kernel, std::atomic<int> (&known)[64][9], int threads, int smem, int cluster) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) { cudaGetLastError(); return kSms / cluster; }
  std::atomic<int>* slot = device < 64 ? &known[device][cluster] : nullptr;
  int n = slot ? slot->load(std::memory_order_relaxed) : 0;
  if (n > 0) return n;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)cluster * 1024);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)cluster;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
      cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    return std::max(1, kSms / cluster);
  }
  if (slot) slot->store(n, std::memory_order_relaxed);
  return n;
}
template <int BN, bool PAIR>
static int wgrad_at_once(int cluster) {
  static std::atomic<int> known[64][9];
  return clusters_at_once(mx_weight_grad_kernel<BN, PAIR>, known, kWgradThreads, WgradSmem<BN, PAIR>::kBytes, cluster);
}

template <int BN, bool PAIR>
static int run_wgrad(const CUtensorMap& codes, const CUtensorMap& grad, const WgradArgs& a, cudaStream_t st) {
  static std::atomic<uint64_t> raised{0};
  const int ctas = PAIR ? 2 : 1;
  return launch_tc(mx_weight_grad_kernel<BN, PAIR>, raised, kWgradThreads, WgradSmem<BN, PAIR>::kBytes, (int64_t)a.k_tiles * a.n_tiles * a.splits * ctas,
                   a.part ? ctas : a.splits * ctas, st, codes, grad, a);
}

// Tile and split of a weight gradient: the fewest nanoseconds, counted as rounds of what runs together times
// (steps times what a step takes with this tile + start and output), and when split either the exchange in a cluster (1.2 us
// and 33 ns to a column of a CTA's share) or the parts' way through memory and the second launch; all measured
// (1024 x 1024 x 1024: 9.8 us unsplit in 128 x 64, 11.9 in 256 x 256 with the sum in three).
struct WgradPlan {
  int bn, ctas, splits;
  bool joined;                            // the parts are joined by join_parts_kernel
  int64_t k_tiles, n_tiles;
};
static WgradPlan plan_wgrad(int64_t tokens, int64_t n, int64_t k, int pieces) {
  const int64_t steps = (tokens + kTok - 1) / kTok * pieces;
  struct Shape { int bn, ctas; double step, fixed; int (*at_once)(int); };
  static const Shape shapes[] = {{512, 2, 560, 6000, wgrad_at_once<512, true>},
                                 {256, 2, 400, 5000, wgrad_at_once<256, true>},
                                 {128, 1, 380, 4500, wgrad_at_once<128, false>},
                                 {64, 1, 360, 4000, wgrad_at_once<64, false>}};
  WgradPlan p{};
  double best = 1e300;
  for (const Shape& c : shapes) {
    const int64_t k_tiles = (k + 128 * c.ctas - 1) / (128 * c.ctas), n_tiles = (n + c.bn - 1) / c.bn, tiles = k_tiles * n_tiles;
    for (int s = 1; s * c.ctas <= 8; ++s) {
      if (s > steps || (s > 1 && c.bn > 256)) continue;      // a split tile has to fit into shared memory
      const int at_once = c.at_once(s * c.ctas);
      const double cost = (double)((tiles + at_once - 1) / at_once) * ((double)((steps + s - 1) / s) * c.step + c.fixed + (s > 1 ? 1200 + 33.0 * c.bn / s : 0));
      if (cost < best) { best = cost; p = {c.bn, c.ctas, s, false, k_tiles, n_tiles}; }
    }
    const int64_t s = std::min<int64_t>(c.at_once(c.ctas) / tiles, steps / 2);
    if (s >= 2 && s * n * k <= ((int64_t)1 << 26)) {
      const double cost = (double)((steps + s - 1) / s) * c.step + c.fixed + 3500 + (double)(s * n * k) * 8 / 8000;     // written and read; fitted to parts that stay in L2
      if (cost < best) { best = cost; p = {c.bn, c.ctas, (int)s, true, k_tiles, n_tiles}; }
    }
  }
  return p;
}

template <int BN>
static int run_fp4(const CUtensorMap& ma, const CUtensorMap& mb, const Fp4Args& a, cudaStream_t st) {
  static std::atomic<uint64_t> raised{0};
  return launch_tc(mx_fp4_kernel<BN>, raised, kFp4Threads, Fp4Smem<BN>::kBytes, (int64_t)a.n_tiles * a.m_tiles * a.splits, a.splits, st, ma, mb, a);
}

template <int BN>
static int fp4_at_once(int cluster) {
  static std::atomic<int> known[64][9];
  return clusters_at_once(mx_fp4_kernel<BN>, known, kFp4Threads, Fp4Smem<BN>::kBytes, cluster);
}
static int fp4_pairs_at_once() {
  static std::atomic<int> known[64][9];
  return clusters_at_once(mx_fp4_pair_kernel, known, kPairThreads, PairSmem::kBytes, 2);
}

// Tile and split of an MXFP4 product, by the microseconds that were measured for each: a start, then rounds of what runs
// together.  Unsplit tiles run two to an SM and slow each other down; clusters run one CTA to an SM.
// (4096 x 4096 x 4096: 45 us in 128 x 128 tiles, 38 in pairs; 2048 x 4096 x 4096: 23 and 25; 1 x 4096 x 4096:
// 8.9 unsplit, 6.4 in four.)
struct Fp4Plan {
  int bm, splits;                         // bm: rows of a to a tile, 384 in pairs
};
static Fp4Plan plan_fp4(int64_t m, int64_t n, int steps) {
  const int64_t n_tiles = (n + 127) / 128;
  const int width = m <= 32 ? 32 : m <= 64 ? 64 : 128;      // narrow ones only for a single tile
  const int64_t tiles = n_tiles * ((m + width - 1) / width);
  Fp4Plan p{width, 1};
  double best = 1e300;
  for (int s = 1; s <= 8 && s <= steps; ++s) {
    const int at_once = s == 1 ? 2 * kSms : width == 128 ? fp4_at_once<128>(s) : width == 64 ? fp4_at_once<64>(s) : fp4_at_once<32>(s);
    const double both = s > 1 ? 0 : std::min(1.0, std::max(0.0, (double)(tiles - kSms) / kSms));     // how far tiles share an SM
    const double round = (double)((steps + s - 1) / s) * (0.34 + 0.15 * both) + (s > 1 ? 3.0 : 1.2 + 1.5 * both);
    const double cost = (s > 1 ? 2.0 : 2.5) + (double)((tiles + at_once - 1) / at_once) * round;
    if (cost < best) { best = cost; p.splits = s; }
  }
  if (m > 128) {
    const int64_t pair_tiles = (n + 255) / 256 * ((m + 383) / 384);
    const int at_once = fp4_pairs_at_once();
    if (3.5 + (double)((pair_tiles + at_once - 1) / at_once) * (steps * 0.5 + 3.0) < best) p = {384, 1};
  }
  return p;
}

static int pieces_of(int dtype) { return dtype == RT_F32 ? 3 : dtype == RT_F16 ? 2 : 1; }
static bool taken_as_is(const void* p, int dtype, int64_t ld) { return dtype == RT_BF16 && aligned16(p, ld, 2); }

}  // namespace rt

using namespace rt;

extern "C" int64_t rt_mx_weight_grad_workspace(const void* grad_out, int grad_dtype, int64_t ld_grad, int64_t tokens, int64_t n, int64_t k) {
  if (!dtype_ok(grad_dtype)) return fail(RT_E_DTYPE, "dtype code must be 0 (bf16), 1 (f32) or 2 (f16)");
  if (int rc = mx_check_shape(tokens, k)) return rc;
  if (int rc = mx_check_shape(tokens, n)) return rc;
  if (tokens == 0 || n == 0 || k == 0) return 0;
  const int pieces = taken_as_is(grad_out, grad_dtype, ld_grad) ? 0 : pieces_of(grad_dtype);
  const WgradPlan plan = plan_wgrad(tokens, n, k, std::max(1, pieces));
  return pad_to(pieces * tokens * pad_to(n, 8) * 2, 16) + (plan.joined ? plan.splits * n * pad_to(k, 4) * 4 : 0);
}

extern "C" int rt_mx_weight_grad_plan(const void* grad_out, int grad_dtype, int64_t ld_grad, int64_t tokens, int64_t n, int64_t k, rt_mx_plan* plan) {
  if (!plan) return fail(RT_E_NULL, "plan must be non-null");
  if (!dtype_ok(grad_dtype)) return fail(RT_E_DTYPE, "dtype code must be 0 (bf16), 1 (f32) or 2 (f16)");
  if (int rc = mx_check_shape(tokens, k)) return rc;
  if (int rc = mx_check_shape(tokens, n)) return rc;
  *plan = rt_mx_plan{};
  if (tokens == 0 || n == 0 || k == 0) return 0;
  const WgradPlan p = plan_wgrad(tokens, n, k, taken_as_is(grad_out, grad_dtype, ld_grad) ? 1 : pieces_of(grad_dtype));
  *plan = {p.bn, p.ctas, p.splits, p.joined};
  return 0;
}

extern "C" int rt_mxfp4_matmul_plan(int64_t m, int64_t n, int64_t k, rt_mx_plan* plan) {
  if (!plan) return fail(RT_E_NULL, "plan must be non-null");
  if (int rc = mx_check_shape(m, k)) return rc;
  if (int rc = mx_check_shape(n, k)) return rc;
  *plan = rt_mx_plan{};
  if (m == 0 || n == 0 || k == 0) return 0;
  const Fp4Plan p = plan_fp4(m, n, (int)((pad_to(k, kMxBlock) + kStepK - 1) / kStepK));
  *plan = {p.bm, p.bm == 384 ? 2 : 1, p.splits, 0};
  return 0;
}

extern "C" int rt_mx_weight_grad(const void* grad_out, int grad_dtype, int64_t ld_grad, const void* codes, const void* scales,
                                 int64_t tokens, int64_t n, int64_t k, void* out, int out_dtype, int64_t ld_out, int accumulate,
                                 void* workspace, int64_t workspace_bytes, void* cuda_stream) {
  if (int rc = mx_check_shape(tokens, k)) return rc;
  if (int rc = mx_check_shape(tokens, n)) return rc;
  if (n == 0 || k == 0) return 0;
  if (int rc = check_out(out, out_dtype, k, ld_out)) return rc;
  if (!dtype_ok(grad_dtype)) return fail(RT_E_DTYPE, "dtype code must be 0 (bf16), 1 (f32) or 2 (f16)");
  cudaStream_t st = (cudaStream_t)cuda_stream;
  if (tokens == 0) {                        // an empty sum
    const size_t size = dtype_size(out_dtype);
    if (!accumulate) RT_CUDA(cudaMemset2DAsync(out, ld_out * size, 0, k * size, n, st));
    return 0;
  }
  if (!grad_out) return fail(RT_E_NULL, "grad_out must be non-null");
  if (ld_grad < n || ld_grad > ((int64_t)1 << 38)) return fail(RT_E_SIZE, "row stride of grad_out must be >= n and at most 2^38");
  if ((uintptr_t)grad_out % dtype_size(grad_dtype)) return fail(RT_E_ALIGN, "grad_out is not aligned to its element size");
  if (int rc = mx_check_codes(codes, scales)) return rc;
  const int64_t need = rt_mx_weight_grad_workspace(grad_out, grad_dtype, ld_grad, tokens, n, k);
  if (need > 0) {
    if (!workspace || workspace_bytes < need) return fail(RT_E_CONFIG, "workspace is smaller than rt_mx_weight_grad_workspace says");
    if ((uintptr_t)workspace & 15) return fail(RT_E_ALIGN, "workspace must be 16-byte aligned");
  }

  const int64_t np = pad_to(n, 8), kp = pad_to(k, kMxBlock);
  const bool spread = !taken_as_is(grad_out, grad_dtype, ld_grad);
  const int pieces = spread ? pieces_of(grad_dtype) : 1;
  const WgradPlan plan = plan_wgrad(tokens, n, k, pieces);
  WgradArgs a{};
  a.scales = (const uint8_t*)scales;
  a.ld_scales = pad_to(kp / kMxBlock, 4);
  a.tokens = (int)tokens;
  a.token_steps = (int)((tokens + kTok - 1) / kTok);
  a.pieces = pieces;
  a.out = {out, ld_out, (int)n, (int)k, out_dtype, accumulate != 0, aligned16(out, ld_out, dtype_size(out_dtype))};

  const OutMatrix result = a.out;
  a.splits = plan.splits;
  a.k_tiles = (int)plan.k_tiles;
  a.n_tiles = (int)plan.n_tiles;
  if (plan.k_tiles * plan.n_tiles * a.splits * plan.ctas > 0x7FFFFFFFll) return fail(RT_E_SIZE, "n * k is too large");
  const int64_t k4 = pad_to(k, 4);
  if (plan.joined) {                        // the parts lie behind the planes
    a.part = n * k4 * 4;
    a.out = {(uint8_t*)workspace + (need - a.splits * a.part), k4, (int)n, (int)k4, RT_F32, 0, 1};
  }

  CUtensorMap map_codes, map_grad;
  {
    const uint64_t dims[2] = {(uint64_t)kp, (uint64_t)tokens}, strides[1] = {(uint64_t)kp};
    const uint32_t box[2] = {128, (uint32_t)kTok};
    if (int rc = make_map(&map_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  }
  {
    const int64_t ld = spread ? np : ld_grad;
    const uint64_t dims[3] = {(uint64_t)n, (uint64_t)tokens, (uint64_t)pieces}, strides[2] = {(uint64_t)ld * 2, (uint64_t)(spread ? tokens * np * 2 : ld * 2)};
    const uint32_t box[3] = {64, (uint32_t)kTok, 1};
    if (int rc = make_map(&map_grad, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, spread ? workspace : grad_out, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  }
  if (spread) {
    if (grad_dtype == RT_F32) run_spread<RT_F32, 3>(grad_out, ld_grad, tokens, n, workspace, st);
    else if (grad_dtype == RT_F16) run_spread<RT_F16, 2>(grad_out, ld_grad, tokens, n, workspace, st);
    else run_spread<RT_BF16, 1>(grad_out, ld_grad, tokens, n, workspace, st);
    if (int rc = launched()) return rc;
  }
  if (int rc = plan.bn == 512   ? run_wgrad<512, true>(map_codes, map_grad, a, st)
               : plan.bn == 256 ? run_wgrad<256, true>(map_codes, map_grad, a, st)
               : plan.bn == 128 ? run_wgrad<128, false>(map_codes, map_grad, a, st)
                                : run_wgrad<64, false>(map_codes, map_grad, a, st))
    return rc;
  if (!plan.joined) return 0;
  const int64_t quads = n * (k4 / 4);
  join_parts_kernel<<<(unsigned)((quads + 255) / 256), 256, 0, st>>>((const float4*)a.out.p, quads, a.splits, FastDiv::of((uint32_t)(k4 / 4)), result);
  return launched();
}

extern "C" int rt_mx_wait_faults(uint32_t* count) {
  if (!count) return fail(RT_E_NULL, "count must be non-null");
  unsigned int v = 0;
  RT_CUDA(cudaMemcpyFromSymbol(&v, g_wait_faults, sizeof v));
  *count = v;
  return 0;
}

extern "C" int rt_mxfp4_matmul(const void* a_codes, const void* a_scales, const void* b_codes, const void* b_scales, int64_t m,
                               int64_t n, int64_t k, void* out, int out_dtype, int64_t ld_out, void* cuda_stream) {
  if (int rc = mx_check_shape(m, k)) return rc;
  if (int rc = mx_check_shape(n, k)) return rc;
  if (m == 0 || n == 0) return 0;
  if (int rc = check_out(out, out_dtype, n, ld_out)) return rc;
  cudaStream_t st = (cudaStream_t)cuda_stream;
  if (k == 0) {                             // an empty sum
    const size_t size = dtype_size(out_dtype);
    RT_CUDA(cudaMemset2DAsync(out, ld_out * size, 0, n * size, m, st));
    return 0;
  }
  if (int rc = mx_check_codes(a_codes, a_scales)) return rc;
  if (int rc = mx_check_codes(b_codes, b_scales)) return rc;
  const int64_t kp = pad_to(k, kMxBlock);
  Fp4Args a{};
  a.a_scales = (const uint8_t*)a_scales;
  a.b_scales = (const uint8_t*)b_scales;
  a.k_padded = (int)kp;
  a.steps = (int)((kp + kStepK - 1) / kStepK);
  a.ktiles = (int)((kp + 127) / 128);
  a.out = {out, ld_out, (int)m, (int)n, out_dtype, 0, aligned16(out, ld_out, dtype_size(out_dtype))};

  const int64_t n_tiles = (n + 127) / 128, pair_tiles = (n + 255) / 256 * ((m + 383) / 384);
  if (pair_tiles > 0x3FFFFFFFll) return fail(RT_E_SIZE, "m * n is too large");
  const auto [bm, splits] = plan_fp4(m, n, a.steps);
  a.splits = splits;
  a.n_tiles = (int)n_tiles;
  a.m_tiles = (int)((m + bm - 1) / bm);
  if (n_tiles * a.m_tiles * splits > 0x7FFFFFFFll) return fail(RT_E_SIZE, "m * n is too large");

  CUtensorMap map_a, map_b;
  const uint64_t strides[1] = {(uint64_t)kp / 2};
  {
    const uint64_t dims[2] = {(uint64_t)kp / 2, (uint64_t)m};
    const uint32_t box[2] = {128, (uint32_t)std::min(bm, 128)};
    if (int rc = make_map(&map_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, a_codes, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  }
  {
    const uint64_t dims[2] = {(uint64_t)kp / 2, (uint64_t)n};
    const uint32_t box[2] = {128, 128};
    if (int rc = make_map(&map_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, b_codes, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  }
  if (bm == 384) {
    CUtensorMap map_a2;
    const uint64_t dims[2] = {(uint64_t)kp / 2, (uint64_t)m};
    const uint32_t box[2] = {128, 64};
    if (int rc = make_map(&map_a2, CU_TENSOR_MAP_DATA_TYPE_UINT8, a_codes, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
    // the scales as rows of tiles, in words: a box is the two tiles of a step, of one or of three row tiles
    CUtensorMap map_sa, map_sb;
    const uint64_t wide[1] = {(uint64_t)a.ktiles * 512};
    const uint64_t dims_a[2] = {(uint64_t)a.ktiles * 128, (uint64_t)(m + 127) / 128}, dims_b[2] = {(uint64_t)a.ktiles * 128, (uint64_t)n_tiles};
    const uint32_t box_a[2] = {256, 3}, box_b[2] = {256, 1};
    if (int rc = make_map(&map_sa, CU_TENSOR_MAP_DATA_TYPE_UINT32, a_scales, 2, dims_a, wide, box_a, CU_TENSOR_MAP_SWIZZLE_NONE)) return rc;
    if (int rc = make_map(&map_sb, CU_TENSOR_MAP_DATA_TYPE_UINT32, b_scales, 2, dims_b, wide, box_b, CU_TENSOR_MAP_SWIZZLE_NONE)) return rc;
    static std::atomic<uint64_t> raised{0};
    a.n_tiles = (int)((n + 255) / 256);
    return launch_tc(mx_fp4_pair_kernel, raised, kPairThreads, PairSmem::kBytes, 2 * std::min<int64_t>(pair_tiles, fp4_pairs_at_once()), 2, st, map_a, map_a2, map_b, map_sa, map_sb, a);
  }
  if (bm == 128) return run_fp4<128>(map_a, map_b, a, st);
  if (bm == 64) return run_fp4<64>(map_a, map_b, a, st);
  return run_fp4<32>(map_a, map_b, a, st);
}
