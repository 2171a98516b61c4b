// The token-policy and 8-bit-activation methods of the CPython module _trl_host (host_policy.cpp), added by host_fast.cpp.
#pragma once
#include <Python.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/jit/frontend/tracer.h>

// Whether torch may be writing down what happens to plain tensors (make_fx, torch.jit.trace): the general path looks closer.
inline bool maybe_recorded() { return c10::impl::TorchDispatchModeTLS::any_modes_set() || torch::jit::tracer::isTracing(); }

extern PyMethodDef trl_policy_methods[];
