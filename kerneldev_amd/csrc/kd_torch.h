// What the C++ routes from torch to the C ABI share: statuses as Python errors,
// and which tensors, modes and cotangents are plain enough for them.
#pragma once
#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <ATen/record_function.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/kdattn.h"

namespace kdt {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

inline PyObject* g_kernel_error = nullptr;  // _lib.KernelError

// A status as the Python layer raises it (_lib.check): ValueError for refused
// arguments, KernelError for the rest
inline void check(int status, const char* what) {
  if (status == KD_OK) return;
  pybind11::gil_scoped_acquire gil;
  std::string msg = std::string(what) + ": " + kd_last_error_string();
  const bool refused = status == KD_ERR_INVALID || status == KD_ERR_UNSUPPORTED;
  if (!refused) msg += " (status " + std::to_string(status) + ")";
  PyErr_SetString(refused ? PyExc_ValueError : g_kernel_error, msg.c_str());
  python_error e;
  e.persist();
  throw e;
}

inline void* stream_on(c10::Device d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }
inline void* stream_of(const Tensor& t) { return stream_on(t.device()); }

// Plain eager tensors: strided GPU tensors with nothing between them and their
// memory (no subclass or mode dispatch, transform, lazy negation or zero, no
// tangent).
inline bool plain(const Tensor& t) {
  using K = c10::DispatchKey;
  static const c10::DispatchKeySet other({K::Python, K::PythonTLSSnapshot, K::Negative, K::Conjugate, K::ZeroTensor,
                                          K::Batched, K::FuncTorchBatched, K::FuncTorchGradWrapper, K::Functionalize});
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.is_nested() &&
         (t.key_set() & other).empty() && !t._fw_grad(0).defined();
}
inline bool plain(const OptTensor& t) { return !t.has_value() || plain(*t); }
inline bool no_dispatch() {  // no dispatch mode, transform or tracer that has to see operations
  using K = c10::DispatchKey;
  return !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
         !c10::impl::tls_is_dispatch_key_included(K::FuncTorchDynamicLayerFrontMode) &&
         !c10::impl::tls_is_dispatch_key_included(K::Functionalize) && !torch::jit::tracer::isTracing();
}
inline bool plain_mode() { return no_dispatch() && at::impl::PythonTorchFunctionTLS::stack_len() == 0; }

// Whether a backward may hand its cotangent to the kernels.  It is whatever the
// nodes behind returned: a batch (is_grads_batched), a tensor with a tangent
// (forward-over-reverse) or a subclass goes through operations that know
// these -- torch's, or the custom op -- and so does everything under a mode that
// was entered for the backward alone.  (Lazy negation and zero tensors are made
// real by the backward itself.)
inline bool plain_cotangent(const Tensor& d) {
  using K = c10::DispatchKey;
  static const c10::DispatchKeySet other({K::Python, K::PythonTLSSnapshot, K::Batched, K::FuncTorchBatched,
                                          K::FuncTorchGradWrapper, K::Functionalize});
  return no_dispatch() && d.is_cuda() && d.layout() == at::kStrided && !d.is_nested() && (d.key_set() & other).empty() &&
         !d._fw_grad(0).defined();
}

// The results of a custom op (attention.py, span_head.py) through the dispatcher
inline variable_list call_op(const char* name, std::vector<c10::IValue> args) {
  const auto op = c10::Dispatcher::singleton().findSchemaOrThrow(name, "");
  op.callBoxed(&args);
  variable_list out;
  for (c10::IValue& r : args) out.push_back(std::move(r).toTensor());
  return out;
}

// Gradients made under create_graph depend on `from` through an op without a
// derivative: going back through them raises, as the custom op does
inline void refuse_second(variable_list& grads, const char* op, const variable_list& from) {
  const auto node = std::make_shared<torch::autograd::Error>(
      std::string("Trying to backward through ") + op + " but no autograd formula was registered.",
      torch::autograd::collect_next_edges(from));
  for (Tensor& g : grads) torch::autograd::set_history(g, node);
}

}  // namespace kdt
