// Host side of the microscaled calls in C++: allocates the results, makes the inputs' device current,
// and calls the C ABI on the current stream.  Shapes, strides and types have been checked by
// ramtorch_b200/microscaling.py, which does the same through ctypes when this module is not built;
// what this saves is Python time (quantize_mxint8 13.0 us a call down to 9.8, weight_grad 16.8 to 10.1, gated_act 36 to 16), which
// is most of a small call.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/extension.h>

#include <vector>

#include "../../include/rt_b200.h"

namespace {

struct Abi {
  decltype(&rt_last_error) last_error = nullptr;
  decltype(&rt_mx_quantize) quantize = nullptr;
  decltype(&rt_mx_dequantize) dequantize = nullptr;
  decltype(&rt_mx_gated_act) gated_act = nullptr;
  decltype(&rt_mx_gated_act_backward) gated_act_backward = nullptr;
  decltype(&rt_mx_weight_grad_workspace) weight_grad_workspace = nullptr;
  decltype(&rt_mx_weight_grad) weight_grad = nullptr;
  decltype(&rt_mxfp4_matmul) matmul = nullptr;
} abi;

template <typename F>
void take(const py::dict& d, const char* name, F& f) {
  f = reinterpret_cast<F>(d[name].cast<uintptr_t>());
}
void init(const py::dict& d) {
  take(d, "rt_last_error", abi.last_error);
  take(d, "rt_mx_quantize", abi.quantize);
  take(d, "rt_mx_dequantize", abi.dequantize);
  take(d, "rt_mx_gated_act", abi.gated_act);
  take(d, "rt_mx_gated_act_backward", abi.gated_act_backward);
  take(d, "rt_mx_weight_grad_workspace", abi.weight_grad_workspace);
  take(d, "rt_mx_weight_grad", abi.weight_grad);
  take(d, "rt_mxfp4_matmul", abi.matmul);
}

void check(int rc, const char* what) {
  if (rc == 0) return;
  const std::string text = std::string(what) + " failed (" + std::to_string(rc) + "): " + abi.last_error();
  if (rc < 0) throw py::value_error(text);
  throw std::runtime_error(text);
}

int code(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? RT_BF16 : t.scalar_type() == at::kFloat ? RT_F32 : RT_F16;
}
at::ScalarType type_of(int dtype) { return dtype == RT_BF16 ? at::kBFloat16 : dtype == RT_F32 ? at::kFloat : at::kHalf; }
at::Tensor empty(at::IntArrayRef size, at::ScalarType type, const c10::Device& device) {
  return at::detail::empty_cuda(size, type, device, std::nullopt);
}
void* stream(const c10::Device& device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }
int64_t pad(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// codes and scales of a matrix, laid out as include/rt_b200.h says
std::pair<at::Tensor, at::Tensor> room(int format, int64_t rows, int64_t cols, const c10::Device& device) {
  const int64_t wide = pad(cols, 32), blocks = wide / 32;
  if (format == RT_MXINT8) return {empty({rows, wide}, at::kChar, device), empty({rows, pad(blocks, 4)}, at::kByte, device)};
  return {empty({rows, wide / 2}, at::kByte, device), empty({pad(rows, 128) / 128, pad(blocks, 4) / 4, 32, 4, 4}, at::kByte, device)};
}

py::tuple quantize(const at::Tensor& x, int64_t rows, int64_t cols, int64_t ld, int format, bool transpose, bool stochastic, uint64_t seed,
                   uint32_t tensor_id, uint32_t step) {
  const c10::cuda::CUDAGuard guard(x.device());
  auto [codes, scales] = room(format, transpose ? cols : rows, transpose ? rows : cols, x.device());
  const rt_mx_draws draws{seed, tensor_id, step};
  check(abi.quantize(x.data_ptr(), code(x), rows, cols, ld, format, transpose, codes.data_ptr(), scales.data_ptr(), stochastic ? &draws : nullptr,
                     stream(x.device())), "rt_mx_quantize");
  return py::make_tuple(codes, scales);
}

at::Tensor dequantize(int format, const at::Tensor& codes, const at::Tensor& scales, int64_t rows, int64_t cols, const std::vector<int64_t>& shape, int dtype) {
  const c10::cuda::CUDAGuard guard(codes.device());
  at::Tensor out = empty(shape, type_of(dtype), codes.device());
  check(abi.dequantize(format, codes.data_ptr(), scales.data_ptr(), rows, cols, out.data_ptr(), dtype, cols, stream(codes.device())), "rt_mx_dequantize");
  return out;
}

py::tuple gated_act(const at::Tensor& gate, int64_t ld_gate, const at::Tensor& up, int64_t ld_up, int64_t rows, int64_t cols, int act) {
  const c10::cuda::CUDAGuard guard(gate.device());
  at::Tensor h = empty(gate.sizes(), gate.scalar_type(), gate.device());
  auto [gc, gs] = room(RT_MXINT8, rows, cols, gate.device());
  auto [uc, us] = room(RT_MXINT8, rows, cols, gate.device());
  check(abi.gated_act(gate.data_ptr(), ld_gate, up.data_ptr(), ld_up, code(gate), rows, cols, act, h.data_ptr(), cols, gc.data_ptr(), gs.data_ptr(),
                      uc.data_ptr(), us.data_ptr(), stream(gate.device())), "rt_mx_gated_act");
  return py::make_tuple(h, gc, gs, uc, us);
}

py::tuple gated_act_backward(const at::Tensor& grad, int64_t ld, int64_t rows, int64_t cols, int act, const at::Tensor& gc, const at::Tensor& gs,
                             const at::Tensor& uc, const at::Tensor& us) {
  const c10::cuda::CUDAGuard guard(grad.device());
  at::Tensor dgate = empty(grad.sizes(), grad.scalar_type(), grad.device()), dup = empty(grad.sizes(), grad.scalar_type(), grad.device());
  check(abi.gated_act_backward(grad.data_ptr(), ld, code(grad), rows, cols, act, gc.data_ptr(), gs.data_ptr(), uc.data_ptr(), us.data_ptr(),
                               dgate.data_ptr(), cols, dup.data_ptr(), cols, stream(grad.device())), "rt_mx_gated_act_backward");
  return py::make_tuple(dgate, dup);
}

at::Tensor weight_grad(const at::Tensor& grad, int64_t ld, const at::Tensor& codes, const at::Tensor& scales, int64_t tokens, int64_t n, int64_t k,
                       const std::optional<at::Tensor>& into, int64_t ld_out, int dtype, bool accumulate) {
  const c10::cuda::CUDAGuard guard(grad.device());
  at::Tensor out = into ? *into : empty({n, k}, type_of(dtype), grad.device());
  const int64_t need = abi.weight_grad_workspace(grad.data_ptr(), code(grad), ld, tokens, n, k);
  if (need < 0) check((int)need, "rt_mx_weight_grad_workspace");
  at::Tensor space;
  if (need > 0) space = empty({need}, at::kByte, grad.device());
  check(abi.weight_grad(grad.data_ptr(), code(grad), ld, codes.data_ptr(), scales.data_ptr(), tokens, n, k, out.data_ptr(), code(out), ld_out, accumulate,
                        need > 0 ? space.data_ptr() : nullptr, need, stream(grad.device())), "rt_mx_weight_grad");
  return out;
}

at::Tensor matmul(const at::Tensor& ac, const at::Tensor& as, const at::Tensor& bc, const at::Tensor& bs, int64_t m, int64_t n, int64_t k,
                  const std::vector<int64_t>& shape, int dtype) {
  const c10::cuda::CUDAGuard guard(ac.device());
  at::Tensor out = empty(shape, type_of(dtype), ac.device());
  check(abi.matmul(ac.data_ptr(), as.data_ptr(), bc.data_ptr(), bs.data_ptr(), m, n, k, out.data_ptr(), dtype, n, stream(ac.device())), "rt_mxfp4_matmul");
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("init", &init);
  m.def("quantize", &quantize);
  m.def("dequantize", &dequantize);
  m.def("gated_act", &gated_act);
  m.def("gated_act_backward", &gated_act_backward);
  m.def("weight_grad", &weight_grad);
  m.def("matmul", &matmul);
}
