// Calls of an operator from Python that do not pass through the dispatcher: Direct<&fn>::call is a CPython function whose `self` is the
// operator's overload in torch.ops.  Plain arguments (dense CUDA tensors of no subclass, int, float, bool, None) go straight to
// fn, which checks them itself; anything else, and a call while a mode, a transform, a tracer or a profiler wants to see operators,
// goes to the overload.  Parsing a call against its schema and boxing it costs as much as the launch (routing of 8 tokens 4.2 us a call, by the
// overload 6.6; 2.5 of both are the launch), and an eager step of one token waits for nothing else.
#pragma once
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/record_function.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <tuple>
#include <utility>

namespace kq_direct {

// keys of a tensor, or of the thread, that somebody else handles before the CUDA kernel
inline bool foreign(c10::DispatchKeySet keys) {
  using K = c10::DispatchKey;
  constexpr c10::DispatchKeySet others({K::Python, K::PythonTLSSnapshot, K::PythonDispatcher, K::Functionalize, K::FuncTorchDynamicLayerFrontMode,
                                        K::FuncTorchDynamicLayerBackMode, K::FuncTorchBatched, K::FuncTorchVmapMode, K::FuncTorchGradWrapper,
                                        K::FuncTorchBatchedDecomposition, K::Batched, K::VmapMode, K::Tracer, K::Conjugate, K::Negative, K::ZeroTensor});
  return keys.has_any(others);
}
inline bool watched() {
  return c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled() || at::hasCallbacks() ||
         foreign(c10::impl::tls_local_dispatch_key_set().included_);
}
inline bool plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.key_set().has(c10::DispatchKey::CUDA) && !foreign(t.key_set());
}

template <typename A> struct Arg;
template <> struct Arg<const at::Tensor&> {
  static bool ok(PyObject* o) { return plain(o); }
  static const at::Tensor& get(PyObject* o) { return THPVariable_Unpack(o); }
};
template <> struct Arg<const std::optional<at::Tensor>&> {
  static bool ok(PyObject* o) { return o == Py_None || plain(o); }
  static std::optional<at::Tensor> get(PyObject* o) { return o == Py_None ? std::nullopt : std::optional<at::Tensor>(THPVariable_Unpack(o)); }
};
template <> struct Arg<int64_t> {
  static bool ok(PyObject* o) {
    int over = 0;
    if (!PyLong_CheckExact(o)) return false;
    PyLong_AsLongLongAndOverflow(o, &over);
    return over == 0;
  }
  static int64_t get(PyObject* o) { return PyLong_AsLongLong(o); }
};
template <> struct Arg<double> {
  static bool ok(PyObject* o) { return PyFloat_CheckExact(o); }
  static double get(PyObject* o) { return PyFloat_AS_DOUBLE(o); }
};
template <> struct Arg<bool> {
  static bool ok(PyObject* o) { return PyBool_Check(o); }
  static bool get(PyObject* o) { return o == Py_True; }
};

inline PyObject* wrap(at::Tensor&& t) { return THPVariable_Wrap(std::move(t)); }      // None where it is not defined
template <typename... T, size_t... I>
PyObject* wrap_all(std::tuple<T...>&& r, std::index_sequence<I...>) {
  PyObject* out = PyTuple_New(sizeof...(T));
  if (!out) return nullptr;
  bool ok = true;
  auto put = [&](size_t i, PyObject* v) {
    ok &= v != nullptr;
    PyTuple_SET_ITEM(out, i, v);
  };
  (put(I, wrap(std::move(std::get<I>(r)))), ...);
  if (!ok) { Py_DECREF(out); return nullptr; }
  return out;
}
template <typename... T> PyObject* wrap(std::tuple<T...>&& r) { return wrap_all(std::move(r), std::index_sequence_for<T...>()); }

template <auto Fn> struct Direct;
template <typename R, typename... A, R (*Fn)(A...)> struct Direct<Fn> {
  template <size_t... I> static PyObject* run(PyObject* self, PyObject* const* args, std::index_sequence<I...>) {
    if (watched() || !(Arg<A>::ok(args[I]) && ...)) return PyObject_Vectorcall(self, args, sizeof...(A), nullptr);
    const std::tuple<decltype(Arg<A>::get(nullptr))...> values(Arg<A>::get(args[I])...);
    std::optional<R> result;
    {
      pybind11::gil_scoped_release others_run;
      result.emplace(std::apply(Fn, values));
    }
    return wrap(std::move(*result));
  }
  static PyObject* call(PyObject* self, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != (Py_ssize_t)sizeof...(A)) return PyObject_Vectorcall(self, args, n, nullptr);
    return run(self, args, std::index_sequence_for<A...>());
    END_HANDLE_TH_ERRORS
  }
};

}  // namespace kq_direct
