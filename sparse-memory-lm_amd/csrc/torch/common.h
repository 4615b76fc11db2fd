// What the wrappers of csrc/torch share: argument checks, streams and workspaces in torch's terms.
#pragma once

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "smlm_pkm.h"

namespace {

using at::Tensor;

inline void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
inline int dtype_of(at::ScalarType t) { return t == at::kFloat ? SMLM_F32 : SMLM_BF16; }
inline bool is_float_type(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }

inline void check(int rc, const char *what) {
  TORCH_CHECK(rc == SMLM_OK, what, " failed with status ", rc, ": ", smlm_pkm_last_error());
}

// t with its values in memory as they are (a view may hold a sign that is yet to be applied).
inline Tensor plain(const Tensor &t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

inline void check_device(const char *name, const Tensor &first, std::initializer_list<const Tensor *> others) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), name, " cannot be traced: a trace would hold its outputs as they were");
  TORCH_CHECK_VALUE(first.is_cuda(), name, ": all tensors must be on a HIP (cuda) device, got ", first.device());
  for (const Tensor *t : others)
    TORCH_CHECK_VALUE(!t->defined() || t->device() == first.device(), name, ": all tensors must be on one device, got ",
                      first.device(), " and ", t->device());
}

inline void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
inline Tensor workspace(const Tensor &like, int64_t bytes) { return at::empty({bytes}, like.options().dtype(at::kByte)); }

}  // namespace
