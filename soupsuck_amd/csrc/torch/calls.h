// What the native entry points share: torch tensors and streams over the C ABI.
#pragma once

#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include "soupsuck_amd.h"

namespace {

using at::Tensor;

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

void check(int rc, const char* name) {
  if (rc == SS_OK) return;
  const std::string text = ss_last_error();
  if (rc == SS_ERR_INVALID_ARGUMENT) TORCH_CHECK_VALUE(false, name, ": ", text);
  TORCH_CHECK(false, name, " failed (", rc, "): ", text);
}

template <class T>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

Tensor empty(at::IntArrayRef sizes, const Tensor& like, at::ScalarType dtype) {
  return at::empty(sizes, like.options().dtype(dtype));
}

Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes ? empty({(int64_t)bytes}, like, at::kByte) : Tensor();
}

}  // namespace
