// Products of microscaled operands: the weight gradient from an 8-bit checkpoint, and the product
// of two MXFP4 matrices.
//
// Simple form: 64 x 64 outputs per CTA, 16 steps of the sum at a time through shared memory, fp32
// multiply-adds in registers.  Every value of either format is exactly an fp32 number, so all that is
// rounded is the sum.
#include <algorithm>

#include "mx_common.cuh"

namespace rt {

int mx_check_shape(int64_t rows, int64_t cols);
int mx_check_codes(const void* codes, const void* scales);

struct FromGradient {       // element (t, i) of a tokens x n gradient
  const void* p;
  int dtype;
  int64_t ld;
  __device__ float operator()(int64_t t, int64_t i) const {
    if (dtype == RT_F32) return static_cast<const float*>(p)[t * ld + i];
    const uint16_t v = static_cast<const uint16_t*>(p)[t * ld + i];
    return dtype == RT_BF16 ? to_f32<RT_BF16>(v) : to_f32<RT_F16>(v);
  }
};
struct FromInt8 {           // element (t, i) of a tokens x k checkpoint
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t ld, ld_scales;
  __device__ float operator()(int64_t t, int64_t i) const {
    return (float)(int8_t)codes[t * ld + i] * scale_of(scales[t * ld_scales + (i >> 5)], 6);
  }
};
struct FromFp4 {            // element (t, i): column t of row i
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t ld;
  int ktiles;
  __device__ float operator()(int64_t t, int64_t i) const {
    const uint32_t c = codes[i * ld + (t >> 1)] >> (4 * (t & 1));
    const float v = __uint_as_float((c & 7u) << 22) * 0x1p126f * scale_of(scales[fp4_scale_at(i, (int)(t >> 5), ktiles)], 0);
    return c & 8u ? -v : v;
  }
};

template <typename A, typename B>
__global__ void __launch_bounds__(256)
simple_product_kernel(const A a, const B b, const int64_t depth, const int64_t rows, const int64_t cols, void* out, const int out_dtype,
                      const int64_t ld, const int accumulate) {
  __shared__ float sa[16][65], sb[16][65];
  const int64_t i0 = (int64_t)blockIdx.y * 64, j0 = (int64_t)blockIdx.x * 64;
  const int ti = threadIdx.x >> 4, tj = threadIdx.x & 15;
  float acc[4][4] = {};
  for (int64_t t0 = 0; t0 < depth; t0 += 16) {
    for (int e = threadIdx.x; e < 1024; e += 256) {
      const int t = e >> 6, i = e & 63;
      const bool live = t0 + t < depth;
      sa[t][i] = live && i0 + i < rows ? a(t0 + t, i0 + i) : 0.f;
      sb[t][i] = live && j0 + i < cols ? b(t0 + t, j0 + i) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 16; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[t][ti + 16 * i], sb[t][tj + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t r = i0 + ti + 16 * i, c = j0 + tj + 16 * j;
      if (r >= rows || c >= cols) continue;
      const int64_t at = r * ld + c;
      if (out_dtype == RT_F32) {
        float* o = static_cast<float*>(out) + at;
        *o = accumulate ? *o + acc[i][j] : acc[i][j];
      } else {
        uint16_t* o = static_cast<uint16_t*>(out) + at;
        if (out_dtype == RT_BF16) *o = of_f32<RT_BF16>(accumulate ? to_f32<RT_BF16>(*o) + acc[i][j] : acc[i][j]);
        else *o = of_f32<RT_F16>(accumulate ? to_f32<RT_F16>(*o) + acc[i][j] : acc[i][j]);
      }
    }
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

}  // namespace rt

using namespace rt;

extern "C" int64_t rt_mx_weight_grad_workspace(const void* grad_out, int grad_dtype, int64_t ld_grad, int64_t tokens, int64_t n, int64_t k) {
  if (!dtype_ok(grad_dtype)) return fail(RT_E_DTYPE, "dtype code must be 0 (bf16), 1 (f32) or 2 (f16)");
  if (int rc = mx_check_shape(tokens, k)) return rc;
  if (int rc = mx_check_shape(tokens, n)) return rc;
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
  if (tokens > 0) {
    if (!grad_out) return fail(RT_E_NULL, "grad_out must be non-null");
    if (ld_grad < n || ld_grad > ((int64_t)1 << 40)) return fail(RT_E_SIZE, "row stride of grad_out must be >= n and at most 2^40");
    if ((uintptr_t)grad_out % dtype_size(grad_dtype)) return fail(RT_E_ALIGN, "grad_out is not aligned to its element size");
    if (int rc = mx_check_codes(codes, scales)) return rc;
  }
  const int64_t kp = pad_to(k, kMxBlock);
  const FromGradient a{grad_out, grad_dtype, ld_grad};
  const FromInt8 b{(const uint8_t*)codes, (const uint8_t*)scales, kp, pad_to(kp / kMxBlock, 4)};
  const dim3 grid((unsigned)((k + 63) / 64), (unsigned)((n + 63) / 64));
  if (grid.y > 65535) return fail(RT_E_SIZE, "n too large");
  simple_product_kernel<<<grid, 256, 0, (cudaStream_t)cuda_stream>>>(a, b, tokens, n, k, out, out_dtype, ld_out, accumulate);
  return launched();
}

extern "C" int rt_mxfp4_matmul(const void* a_codes, const void* a_scales, const void* b_codes, const void* b_scales, int64_t m,
                               int64_t n, int64_t k, void* out, int out_dtype, int64_t ld_out, void* cuda_stream) {
  if (int rc = mx_check_shape(m, k)) return rc;
  if (int rc = mx_check_shape(n, k)) return rc;
  if (m == 0 || n == 0) return 0;
  if (int rc = check_out(out, out_dtype, n, ld_out)) return rc;
  if (k > 0) {
    if (int rc = mx_check_codes(a_codes, a_scales)) return rc;
    if (int rc = mx_check_codes(b_codes, b_scales)) return rc;
  }
  const int64_t kp = pad_to(k, kMxBlock);
  const int kt = (int)((kp + 127) / 128);
  const FromFp4 a{(const uint8_t*)a_codes, (const uint8_t*)a_scales, kp / 2, kt}, b{(const uint8_t*)b_codes, (const uint8_t*)b_scales, kp / 2, kt};
  const dim3 grid((unsigned)((n + 63) / 64), (unsigned)((m + 63) / 64));
  if (grid.y > 65535) return fail(RT_E_SIZE, "m too large");
  simple_product_kernel<<<grid, 256, 0, (cudaStream_t)cuda_stream>>>(a, b, k, m, n, out, out_dtype, ld_out, 0);
  return launched();
}
